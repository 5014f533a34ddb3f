"""The quantised cache and its attention on the device against numpy.

Codes, scales and rotated rows follow from their definitions bit by bit.
Attention is compared with float64 on the same cached values, at 1e-5 of the
largest output. The kernels keep fp32 accuracy: a score is head_dim products
of 22-bit factors or better, summed in fp32, so its error is about 2^-24 of
the root of the sum's squared partial sums (scale * sqrt(128) * 2^-24 * ~8
for N(0, 1) queries and keys: 5e-7), and a relative error of that size in
every weight moves an output by the same part of sqrt(sum w^2) |v|, which is
the size of the outputs themselves; the value sums add 2^-24 sqrt(n) / 2 of
it at n equally weighted positions (3e-6 at 10^4). 1e-5 leaves a factor of
three over the largest of a few thousand outputs.
"""
import math

import numpy as np
import pytest

import attn_ref as ref
from hako_amd.gpu import KV_F16, KV_Q8, HakoGpuError, Rope

pytestmark = pytest.mark.gpu

TUNE_ATTN_PROMPT = 21

TOL = 1e-5
KINDS = [KV_Q8, KV_F16]


def close(got, want, tol=TOL):
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    top = np.nanmax(np.abs(want)) if want.size and not np.isnan(want).all() else 0.0
    err = np.nanmax(np.abs(got - want)) if want.size and not np.isnan(want).all() else 0.0
    assert err <= tol * top, f"error {err:.3g} of {top:.3g}"


def i32(gpu, v):
    return gpu.upload(np.asarray(v, np.int32))


# ── append and read ──

def special_rows(x):
    """Rows that a quantiser meets seldom: zeros, one value, subnormals, huge and tiny ones, ties."""
    hd = x.shape[-1]
    flat = x.reshape(-1, hd)
    flat[0] = 0
    if len(flat) > 8:
        flat[1] = 0
        flat[1, 3] = -5.0
        flat[2] = 1e-40
        flat[3] *= 1e30
        flat[4] *= 1e-30
        flat[5] = np.arange(hd) - hd / 2 + 0.5          # halves: 127 / max is no power of two
        flat[6] = np.where(np.arange(hd) % 2, 127.0, 2.5)   # products that tie
        flat[7] = 2e-38
        flat[8, 7] = 3e38
    return x


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,kvh,H,n,rot,inter,pad", [
    (128, 2, 16, 1, 128, 0, 0), (128, 4, 28, 5, 128, 1, 4), (64, 2, 14, 67, 64, 0, 0), (64, 1, 1, 3, 8, 1, 12),
    (128, 1, 3, 33, 96, 0, 0), (128, 3, 6, 17, 96, 1, 8), (64, 8, 8, 130, 48, 0, 0), (128, 2, 0, 9, 0, 0, 0),
    (64, 5, 10, 2, 32, 1, 0)])
def test_append_and_read(gpu, kind, hd, kvh, H, n, rot, inter, pad):
    rng = np.random.default_rng(hd * n + rot)
    slots, max_seq = 3, 200
    c = ref.Cache(gpu, kind, slots, max_seq, kvh, hd, fill=9)
    D, KV = H * hd, kvh * hd
    ld = D + 2 * KV + pad
    x = rng.standard_normal((n, ld)).astype(np.float32)
    x[:, D + KV:D + 2 * KV] = special_rows(x[:, D + KV:D + 2 * KV].reshape(n, kvh, hd).copy()).reshape(n, KV)
    where = rng.permutation(slots * max_seq)[:n]
    slot, pos = (where // max_seq).astype(np.int32), (where % max_seq).astype(np.int32)
    tab = ref.table(max_seq, rot, stretch=2.0) if rot else None
    dx, ds, dp = gpu.upload(x), i32(gpu, slot), i32(gpu, pos)
    dq = gpu.upload(np.full((n, D + 4), 7, np.float32)) if H else None
    dt = gpu.upload(tab) if rot else None
    gpu.kv_append(c.kv, ds, dp, n, dx.offset(4 * D), dx.offset(4 * (D + KV)), ld,
                  Rope(dt.ptr, max_seq, rot, inter) if rot else None, dx if H else None, dq, H, ld, D + 4)
    k, v = x[:, D:D + KV].reshape(n, kvh, hd), x[:, D + KV:D + 2 * KV].reshape(n, kvh, hd)
    if rot:
        k = ref.rotate(k, tab[pos], rot, inter)
    if H:
        got = gpu.download(dq, np.float32, (n, D + 4))
        np.testing.assert_array_equal(got[:, :D].reshape(n, H, hd), ref.rotate(x[:, :D].reshape(n, H, hd), tab[pos], rot, inter))
        assert (got[:, D:] == 7).all()
    c.k[slot, :, pos], c.ks[slot, :, pos] = ref.rows(k, kind)
    c.v[slot, :, pos], c.vs[slot, :, pos] = ref.rows(v, kind)
    for got, want in zip(c.pull(), (c.k, c.v, c.ks, c.vs)):
        np.testing.assert_array_equal(got, want)   # the rows written and the rows left alone
    # read back, some tokens outside the cache
    pos[n // 2] = max_seq if n > 1 else pos[0]
    dp2, dk, dv = i32(gpu, pos), *(gpu.upload(np.full((n, KV + pad), 3, np.float32)) for _ in range(2))
    gpu.kv_read(c.kv, ds, dp2, n, dk, dv, KV + pad)
    for buf, codes, scales in ((dk, c.k, c.ks), (dv, c.v, c.vs)):
        want = np.full((n, KV + pad), 3, np.float32)
        for i in range(n):
            if pos[i] < max_seq:
                want[i, :KV] = (codes[slot[i], :, pos[i]].astype(np.float32) * scales[slot[i], :, pos[i], None]).reshape(-1)
        np.testing.assert_array_equal(gpu.download(buf, np.float32, want.shape), want)
    for b in (dx, ds, dp, dp2, dq, dt, dk, dv):
        if b:
            b.free()
    c.free()


@pytest.mark.parametrize("kind", KINDS)
def test_append_leaves_out_and_in_place(gpu, kind):
    """Padding (-1), slots and positions past the cache or the table: nothing of the token is written."""
    hd, kvh, H, n, max_seq = 128, 2, 4, 9, 64
    rng = np.random.default_rng(3)
    c = ref.Cache(gpu, kind, 2, max_seq, kvh, hd, fill=5)
    KV, D = kvh * hd, H * hd
    q, k, v = (rng.standard_normal((n, w)).astype(np.float32) for w in (D, KV, KV))
    slot = np.array([0, -1, 1, 2, 0, 1, 2 ** 31 - 1, 1, 0], np.int32)
    pos = np.array([0, 1, -1, 3, 63, 64, 5, 50, -2 ** 31], np.int32)
    tab = ref.table(48, hd)
    ok = [0]   # 63 and 50 lie past the table's 48 positions
    bufs = [gpu.upload(a) for a in (q, k, v, slot, pos, tab)]
    dq, dk, dv, ds, dp, dt = bufs
    gpu.kv_append(c.kv, ds, dp, n, dk, dv, KV, Rope(dt.ptr, 48, hd, 0), dq, dq, H, D, D)
    want = q.copy()
    want[ok] = ref.rotate(q[ok].reshape(-1, H, hd), tab[pos[ok]], hd, 0).reshape(-1, D)
    np.testing.assert_array_equal(gpu.download(dq, np.float32, q.shape), want)
    kk = ref.rotate(k[ok].reshape(-1, kvh, hd), tab[pos[ok]], hd, 0)
    c.k[slot[ok], :, pos[ok]], c.ks[slot[ok], :, pos[ok]] = ref.rows(kk, kind)
    c.v[slot[ok], :, pos[ok]], c.vs[slot[ok], :, pos[ok]] = ref.rows(v[ok].reshape(-1, kvh, hd), kind)
    for got, w in zip(c.pull(), (c.k, c.v, c.ks, c.vs)):
        np.testing.assert_array_equal(got, w)
    for b in bufs:
        b.free()
    c.free()


@pytest.mark.parametrize("kind", KINDS)
def test_rows_that_are_not_finite(gpu, kind):
    hd, max_seq = 64, 8
    c = ref.Cache(gpu, kind, 1, max_seq, 1, hd, fill=0)
    x = np.random.default_rng(0).standard_normal((4, hd)).astype(np.float32)
    x[0, 5], x[1, 63], x[2, 0] = np.nan, np.inf, -np.inf
    d, p, s = gpu.upload(x), i32(gpu, range(4)), i32(gpu, [0] * 4)
    gpu.kv_append(c.kv, s, p, 4, d, d, hd)
    k, _, ks, _ = c.pull()
    assert np.isnan(ks[0, 0, :3]).all() and (k[0, 0, :3] == 0).all() and np.isfinite(ks[0, 0, 3])
    out = gpu.alloc(x.nbytes)
    gpu.kv_read(c.kv, s, p, 4, out, None, hd)
    got = gpu.download(out, np.float32, x.shape)
    assert np.isnan(got[:3]).all() and np.isfinite(got[3]).all()
    # a token that sees such a row answers NaN, one that does not is untouched by it
    c.k[:], c.v[:], c.ks[:], c.vs[:] = c.pull()
    q, ln, o = gpu.upload(x[3]), i32(gpu, [4]), gpu.alloc(4 * hd)
    gpu.attn_decode(o, hd, q, hd, c.kv, s, ln, 1, 1, 0.125)
    assert np.isnan(gpu.download(o, np.float32, (hd,))).all()
    for b in (d, p, s, out, q, ln, o):
        b.free()
    c.free()


# ── attention of single tokens ──

def run_decode(gpu, c, q, slot, lens, scale, ps=0, pl=0, pad=0, in_place=False):
    n, H, hd = q.shape
    ld = H * hd + pad
    host = np.full((n, ld), 3, np.float32)
    host[:, :H * hd] = q.reshape(n, -1)
    dq = gpu.upload(host)
    do = dq if in_place else gpu.upload(np.full((n, H * hd + 8), 11, np.float32))
    ldo = ld if in_place else H * hd + 8
    ds, dl = None if slot is None else i32(gpu, slot), i32(gpu, lens)
    gpu.attn_decode(do, ldo, dq, ld, c.kv, ds, dl, n, H, scale, ps, pl)
    got = gpu.download(do, np.float32, (n, ldo))
    assert (got[:, H * hd:] == (3 if in_place else 11)).all()
    for b in {dq, do, dl} | ({ds} if ds else set()):
        b.free()
    return got[:, :H * hd].reshape(n, H, hd)


def want_decode(c, q, slot, lens, scale, ps=0, pl=0):
    K, V = c.values()
    out = []
    for i, m in enumerate(lens):
        s = i if slot is None else slot[i]
        m = min(max(m, 0), c.max_seq) if 0 <= s < c.slots else 0
        out.append(ref.attend(q[i], K, V, s, m, scale, ps, pl))
    return np.stack(out)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,kvh,G,max_seq,lens", [
    (128, 2, 8, 1100, [1025]), (128, 4, 7, 700, [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 700, 0]),
    (64, 2, 7, 333, [333, 0, 332, 5]), (64, 1, 1, 64, [64, 1]), (128, 1, 16, 300, [299, 64, 300]),
    (128, 8, 1, 257, [257, 256, 255]), (64, 3, 5, 1, [1, 0]), (128, 2, 3, 5000, [5000, 4097]),
    (64, 4, 16, 2100, [2100, 1999, 3]), (128, 1, 1, 20000, [19999])])
def test_decode(gpu, kind, hd, kvh, G, max_seq, lens):
    rng = np.random.default_rng(max_seq + G)
    c = ref.Cache(gpu, kind, len(lens), max_seq, kvh, hd, rng)
    q = rng.standard_normal((len(lens), kvh * G, hd)).astype(np.float32)
    scale = 1 / math.sqrt(hd)
    close(run_decode(gpu, c, q, None, lens, scale), want_decode(c, q, None, lens, scale))
    c.free()


@pytest.mark.parametrize("kind", KINDS)
def test_decode_slots_strides_in_place(gpu, kind):
    """Slots in any order, one twice, one outside; lengths past the cache and below 0."""
    rng = np.random.default_rng(8)
    c = ref.Cache(gpu, kind, 5, 150, 2, 128, rng)
    slot = [4, 0, 4, 5, -1, 2, 1, 2 ** 31 - 1]
    lens = [150, 77, 3, 20, 20, 2 ** 31 - 1, -5, 9]
    q = rng.standard_normal((len(slot), 12, 128)).astype(np.float32)
    want = want_decode(c, q, slot, lens, 0.07)
    assert (want[[3, 4, 6, 7]] == 0).all()
    close(run_decode(gpu, c, q, slot, lens, 0.07, pad=20), want)
    close(run_decode(gpu, c, q, slot, lens, 0.07, pad=4, in_place=True), want)
    c.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,kvh,G,n,pl,own", [
    (128, 4, 7, 9, 130, 70), (64, 2, 4, 3, 64, 1), (128, 2, 8, 16, 1000, 33), (128, 1, 16, 2, 1, 200),
    (64, 1, 1, 40, 517, 0), (128, 2, 3, 1, 300, 20), (128, 1, 5, 67, 64, 64), (64, 2, 16, 20, 2049, 5)])
def test_decode_prefix(gpu, kind, hd, kvh, G, n, pl, own):
    """A prefix in one slot; some sequences end inside it, one sees nothing."""
    rng = np.random.default_rng(pl)
    max_seq = pl + own + 40
    c = ref.Cache(gpu, kind, n + 1, max_seq, kvh, hd, rng)
    lens = [pl + 1 + (i * 7) % (own + 1) for i in range(n)]
    if n > 2:
        lens[1], lens[2] = pl // 2, 0
    q = rng.standard_normal((n, kvh * G, hd)).astype(np.float32)
    want = want_decode(c, q, None, lens, 0.1, n, pl)
    close(run_decode(gpu, c, q, None, lens, 0.1, n, pl), want)
    # the sequences' own rows below the prefix are not read
    c.k[:n, :, :pl], c.v[:n, :, :pl], c.ks[:n, :, :pl], c.vs[:n, :, :pl] = 1, 1, np.nan, np.nan
    c.push()
    close(run_decode(gpu, c, q, None, lens, 0.1, n, pl), want)
    c.free()


@pytest.mark.parametrize("kind", KINDS)
def test_decode_does_not_read_past_the_end(gpu, kind):
    """Rows past a length may hold anything: NaN scales, and NaN and infinite halves."""
    rng = np.random.default_rng(2)
    c = ref.Cache(gpu, kind, 3, 400, 2, 128, rng)
    lens = [37, 0, 390]
    q = rng.standard_normal((3, 8, 128)).astype(np.float32)
    want = want_decode(c, q, None, lens, 0.09)
    for i, m in enumerate(lens):
        c.ks[i, :, m:], c.vs[i, :, m:] = np.nan, np.inf
        c.k[i, :, m:], c.v[i, :, m:] = (127, -127) if kind == KV_Q8 else (np.nan, np.inf)
    c.push()
    close(run_decode(gpu, c, q, None, lens, 0.09), want)
    c.free()


def test_decode_large_scores(gpu):
    """Scores of several hundred: the weights are those of the largest, with no overflow; and a flat row."""
    rng = np.random.default_rng(12)
    c = ref.Cache(gpu, KV_Q8, 2, 300, 1, 64, rng)
    q = np.stack([rng.standard_normal((2, 64)) * 300, np.zeros((2, 64))]).astype(np.float32)
    want = want_decode(c, q, None, [300, 300], 0.125)
    got = run_decode(gpu, c, q, None, [300, 300], 0.125)
    # scores of about 300 * 0.125 * 8 = 300 with 2^-23 of error each way: weights off by 300 * 2^-22
    close(got[0], want[0], 300 * 2.0 ** -21)
    close(got[1], want[1])
    c.free()


def test_decode_past_4_gib(gpu):
    """The last slot of a cache of 4.7 GB per array: offsets past 32 bits."""
    import ctypes as C

    from hako_amd.gpu import Kv
    hd, kvh, max_seq, slots, n = 128, 8, 65536, 70, 40
    kv = Kv(KV_Q8, slots, max_seq, kvh, hd)
    codes, scales = gpu.kv_bytes(kv)
    assert codes > 1 << 32
    bufs = [gpu.alloc(b) for b in (codes, codes, scales, scales)]
    kv.k, kv.v, kv.k_scale, kv.v_scale = (b.ptr for b in bufs)
    rng = np.random.default_rng(1)
    x = rng.standard_normal((n, 2, kvh, hd)).astype(np.float32)
    dx, ds, dp = gpu.upload(x), i32(gpu, [slots - 1] * n), i32(gpu, range(n))
    gpu.kv_append(kv, ds, dp, n, dx, dx.offset(4 * kvh * hd), 2 * kvh * hd)
    q = rng.standard_normal((1, 2 * kvh, hd)).astype(np.float32)
    dq, dl, do = gpu.upload(q), i32(gpu, [n]), gpu.alloc(q.nbytes)
    s1 = i32(gpu, [slots - 1])
    gpu.attn_decode(do, q[0].size, dq, q[0].size, kv, s1, dl, 1, 2 * kvh, 0.1)
    ck, cks = ref.rows(x[:, 0], KV_Q8)
    cv, cvs = ref.rows(x[:, 1], KV_Q8)
    K, V = ((a.astype(np.float64) * b.astype(np.float64)[..., None]).transpose(1, 0, 2)[None] for a, b in ((ck, cks), (cv, cvs)))
    want = ref.attend(q[0], K, V, 0, n, 0.1)
    close(gpu.download(do, np.float32, want.shape), want)
    h = [np.array([v], np.int32) for v in (slots - 1, n - 1, 1)]
    gpu.attn_prompt(do, q[0].size, dq, q[0].size, kv, *h, 1, 2 * kvh, 0.1)
    close(gpu.download(do, np.float32, want.shape), want)
    for b in bufs + [dx, ds, dp, dq, dl, do, s1]:
        b.free()


# ── attention of whole prompts ──

@pytest.fixture(params=[0, 1, 2], ids=["by shape", "direct", "tiled"])
def prompt_kernel(gpu, request):
    gpu.tune(TUNE_ATTN_PROMPT, request.param)
    yield request.param
    gpu.tune(TUNE_ATTN_PROMPT, 0)


def run_prompt(gpu, c, q, slot, start, lens, scale, ps=0, pl=0, pad=0, in_place=False):
    n, H, hd = q.shape
    ld = H * hd + pad
    host = np.full((max(n, 1) + 1, ld), 3, np.float32)
    host[:n, :H * hd] = q.reshape(n, -1)
    dq = gpu.upload(host)
    do = dq if in_place else gpu.upload(np.full(host.shape, 11, np.float32))
    arrays = [None if a is None else np.asarray(a, np.int32) for a in (slot, start, lens)]
    gpu.attn_prompt(do, ld, dq, ld, c.kv, *arrays, len(lens), H, scale, ps, pl)
    got = gpu.download(do, np.float32, host.shape)
    fill = 3 if in_place else 11
    assert (got[n:] == fill).all() and (got[:n, H * hd:] == fill).all()   # the row behind the last, the padding
    for b in {dq, do}:
        b.free()
    return got[:n, :H * hd].reshape(n, H, hd)


def want_prompt(c, q, slot, start, lens, scale, ps=0, pl=0):
    K, V = c.values()
    out, row = [], 0
    for s, (a, m) in enumerate(zip(start, lens)):
        for i in range(m):
            out.append(ref.attend(q[row + i], K, V, s if slot is None else slot[s], a + i + 1, scale, ps, pl))
        row += m
    return np.stack(out)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,kvh,G,max_seq,start,lens", [
    (128, 2, 8, 80, [0], [77]), (128, 4, 7, 600, [0, 200, 0, 63, 64, 65], [130, 77, 0, 1, 65, 17]),
    (64, 2, 7, 300, [0, 31], [257, 129]), (64, 1, 1, 200, [0, 100, 199], [200, 33, 1]), (128, 1, 16, 100, [1], [99]),
    (128, 3, 5, 520, [511, 0], [9, 1]), (64, 8, 2, 128, [0, 0, 0], [128, 127, 1]), (128, 1, 3, 1500, [0], [700]),
    (128, 2, 1, 3000, [2900, 0], [64, 40]), (64, 1, 16, 4200, [4096, 0], [100, 3])])
def test_prompt(gpu, prompt_kernel, kind, hd, kvh, G, max_seq, start, lens):
    rng = np.random.default_rng(max_seq + hd)
    c = ref.Cache(gpu, kind, len(lens), max_seq, kvh, hd, rng)
    q = rng.standard_normal((sum(lens), kvh * G, hd)).astype(np.float32)
    scale = 1 / math.sqrt(hd)
    close(run_prompt(gpu, c, q, None, start, lens, scale), want_prompt(c, q, None, start, lens, scale))
    c.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pl", [1, 63, 64, 100, 190])
def test_prompt_prefix_slots_strides(gpu, prompt_kernel, kind, pl):
    """A prefix in common of any length, a slot named twice, prompts that begin inside the prefix."""
    rng = np.random.default_rng(pl)
    c = ref.Cache(gpu, kind, 4, 400, 2, 128, rng)
    slot, start, lens = [2, 0, 2, 1], [pl, pl + 70, 0, pl // 2], [70, 33, 250, 100]
    q = rng.standard_normal((sum(lens), 6, 128)).astype(np.float32)
    want = want_prompt(c, q, slot, start, lens, 0.08, 3, pl)
    close(run_prompt(gpu, c, q, slot, start, lens, 0.08, 3, pl, pad=12), want)
    close(run_prompt(gpu, c, q, slot, start, lens, 0.08, 3, pl, in_place=True), want)
    c.free()


@pytest.mark.parametrize("kind", KINDS)
def test_prompt_masked_rows(gpu, prompt_kernel, kind):
    """What a token may not see may hold anything: rows past the prompt's end NaN, and a later token's row not finite."""
    rng = np.random.default_rng(5)
    c = ref.Cache(gpu, kind, 2, 200, 1, 128, rng)
    start, lens = [0, 30], [100, 71]
    q = rng.standard_normal((171, 4, 128)).astype(np.float32)
    want = want_prompt(c, q, None, start, lens, 0.09)
    for i in range(2):
        e = start[i] + lens[i]
        c.ks[i, :, e:], c.vs[i, :, e:] = np.nan, np.inf
        c.k[i, :, e:], c.v[i, :, e:] = (127, -127) if kind == KV_Q8 else (np.nan, np.inf)
    c.k[0, :, 90], c.ks[0, :, 90] = 0, np.nan      # as an appended row with a NaN: seen from position 90 on
    c.v[0, :, 70], c.vs[0, :, 70] = 0, np.nan
    want[70:100] = np.nan
    c.push()
    close(run_prompt(gpu, c, q, None, start, lens, 0.09), want)
    c.free()


@pytest.mark.parametrize("kind", KINDS)
def test_prompt_later_rows_do_not_count(gpu, prompt_kernel, kind):
    """A token's output does not depend on the rows after it by a bit, whatever their size."""
    rng = np.random.default_rng(6)
    c = ref.Cache(gpu, kind, 2, 200, 1, 128, rng)
    start, lens, at = [0, 30], [100, 71], 60
    q = rng.standard_normal((171, 4, 128)).astype(np.float32)
    before = [i for i in range(171) if (i if i < 100 else i - 70) < at]
    first = run_prompt(gpu, c, q, None, start, lens, 0.09)
    close(first, want_prompt(c, q, None, start, lens, 0.09))
    c.ks[:, :, at:] *= 2.0 ** 20
    c.vs[:, :, at:] *= 2.0 ** 70
    c.push()
    got = run_prompt(gpu, c, q, None, start, lens, 0.09)
    assert np.isfinite(got).all()
    np.testing.assert_array_equal(got[before], first[before])
    c.free()


@pytest.mark.parametrize("kind", KINDS)
def test_decode_prefix_rows_past_a_length_do_not_count(gpu, kind):
    rng = np.random.default_rng(7)
    c = ref.Cache(gpu, kind, 4, 400, 1, 128, rng)
    lens, pl = [100, 77, 33], 300
    q = rng.standard_normal((3, 4, 128)).astype(np.float32)
    first = run_decode(gpu, c, q, None, lens, 0.09, 3, pl)
    close(first, want_decode(c, q, None, lens, 0.09, 3, pl))
    c.ks[3, :, 100:] *= 2.0 ** 20
    c.vs[3, :, 100:] *= 2.0 ** 70
    c.push()
    np.testing.assert_array_equal(run_decode(gpu, c, q, None, lens, 0.09, 3, pl), first)
    c.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [2.0 ** 70, 2.0 ** -70])
def test_values_of_any_size(gpu, prompt_kernel, kind, size):
    """Large and small values, after rows of zeros and rows that are far smaller."""
    rng = np.random.default_rng(17)
    c = ref.Cache(gpu, kind, 1, 500, 2, 64, rng)
    c.vs *= np.float32(size)
    c.vs[:, :, :70] *= np.float32(2.0 ** -9)
    c.v[:, :, :40], c.vs[:, :, :40] = 0, ref.rows(np.zeros(64, np.float32), kind)[1]
    c.push()
    q = rng.standard_normal((90, 6, 64)).astype(np.float32)
    for start in (0, 45, 410):
        close(run_prompt(gpu, c, q, None, [start], [90], 0.125), want_prompt(c, q, None, [start], [90], 0.125))
    for n in (40, 60, 500):
        close(run_decode(gpu, c, q[:1], None, [n], 0.125), want_decode(c, q[:1], None, [n], 0.125))
    c.free()


def test_prompt_many_sequences(gpu, prompt_kernel):
    """More sequences than one launch takes, most of them short or empty."""
    rng = np.random.default_rng(9)
    n = 300
    c = ref.Cache(gpu, KV_Q8, 40, 30, 1, 64, rng)
    lens = [(i * 5) % 7 if i % 3 else 0 for i in range(n)]
    start, slot = [i % 20 for i in range(n)], [(i * 11) % 40 for i in range(n)]
    q = rng.standard_normal((sum(lens), 2, 64)).astype(np.float32)
    close(run_prompt(gpu, c, q, slot, start, lens, 0.125), want_prompt(c, q, slot, start, lens, 0.125))
    gpu.attn_prompt(*_dummy(gpu, c), c.kv, None, *(np.zeros(2, np.int32) for _ in range(2)), 2, 2, 0.1)   # nothing to do
    gpu.attn_prompt(*_dummy(gpu, c), c.kv, None, None, None, 0, 2, 0.1)
    c.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,kvh,G,start,lens,prefix", [
    (128, 4, 7, [0, 500], [4500, 700], 0),        # whole tiles and parts, in order of length
    (64, 1, 16, [0], [8100], 0),                  # more items than the order's table holds
    (128, 8, 4, [1000, 1000, 1000], [1500, 40, 900], 1000)])
def test_prompt_long(gpu, prompt_kernel, kind, hd, kvh, G, start, lens, prefix):
    """Long prompts, a sample of their tokens against float64: the first, the last, those at tile and chunk borders."""
    if prompt_kernel == 1 and sum(lens) > 5000:
        pytest.skip("the tiled kernel's range")
    rng = np.random.default_rng(hd + G)
    n_seq = len(lens)
    c = ref.Cache(gpu, kind, n_seq + 1, max(a + m for a, m in zip(start, lens)), kvh, hd, rng)
    q = rng.standard_normal((sum(lens), kvh * G, hd)).astype(np.float32)
    got = run_prompt(gpu, c, q, None, start, lens, 1 / math.sqrt(hd), n_seq, prefix)
    assert np.isfinite(got).all()
    K, V = c.values()
    row, at, want = 0, [], []
    for s, (a, m) in enumerate(zip(start, lens)):
        T = 256 // G
        for i in {0, m - 1, m // 2, min(T, m) - 1, min(T, m - 1), max(0, m // T * T - 1), max(0, 64 - a - 1) % m, *rng.integers(0, m, 12)}:
            at.append(row + int(i))
            want.append(ref.attend(q[row + i], K, V, s, a + int(i) + 1, 1 / math.sqrt(hd), n_seq, prefix))
        row += m
    close(got[at], np.stack(want))
    c.free()


def test_decode_many_sequences(gpu):
    """More sequences than CUs, one part each; with and without a prefix."""
    rng = np.random.default_rng(50)
    n = 300
    c = ref.Cache(gpu, KV_Q8, 61, 260, 2, 64, rng)
    slot, lens = [i % 60 for i in range(n)], [(i * 37) % 261 for i in range(n)]
    q = rng.standard_normal((n, 6, 64)).astype(np.float32)
    close(run_decode(gpu, c, q, slot, lens, 0.125), want_decode(c, q, slot, lens, 0.125))
    close(run_decode(gpu, c, q, slot, lens, 0.125, 60, 111), want_decode(c, q, slot, lens, 0.125, 60, 111))
    c.free()


@pytest.mark.parametrize("kind", KINDS)
def test_decode_long_ones_among_many(gpu, kind):
    """Sequences enough for every CU: the long ones in parts, the short ones written at once, in place too."""
    rng = np.random.default_rng(51)
    n = 260
    c = ref.Cache(gpu, kind, 5, 4200, 1, 64, rng)
    slot = [i % 5 for i in range(n)]
    lens = [{3: 4200, 50: 2048, 51: 2049, 100: 0, 101: 4097}.get(i, 1 + (i * 53) % 300) for i in range(n)]
    q = rng.standard_normal((n, 3, 64)).astype(np.float32)
    want = want_decode(c, q, slot, lens, 0.125)
    close(run_decode(gpu, c, q, slot, lens, 0.125), want)
    close(run_decode(gpu, c, q, slot, lens, 0.125, in_place=True), want)
    close(run_decode(gpu, c, q, slot, lens, 0.125, 4, 90), want_decode(c, q, slot, lens, 0.125, 4, 90))
    c.free()


@pytest.mark.parametrize("kind", KINDS)
def test_captured_prompt(gpu, prompt_kernel, kind):
    """An append and a prompt in parts, captured: each replay equals the eager calls on the same rows."""
    hd, kvh, H, n, at = 128, 2, 14, 90, 900
    D, KV = H * hd, kvh * hd
    ld = D + 2 * KV
    rng = np.random.default_rng(60)
    c = ref.Cache(gpu, kind, 2, 1000, kvh, hd, rng)
    tab = ref.table(1000, hd)
    bufs = [gpu.alloc(4 * n * ld), i32(gpu, [1] * n), i32(gpu, range(at, at + n)), gpu.alloc(4 * n * D), gpu.upload(tab)]
    dx, ds, dp, dq, dt = bufs
    host = [np.array([v], np.int32) for v in (1, at, n)]

    def calls():
        gpu.kv_append(c.kv, ds, dp, n, dx.offset(4 * D), dx.offset(4 * (D + KV)), ld, Rope(dt.ptr, 1000, hd, 1), dx, dq, H, ld, D)
        gpu.attn_prompt(dq, D, dq, D, c.kv, *host, 1, H, 0.09)

    gpu.h2d(dx, np.zeros((n, ld), np.float32))
    calls()
    gpu.capture_begin()
    calls()
    graph = gpu.capture_end()
    for _ in range(3):
        y = rng.standard_normal((n, ld)).astype(np.float32)
        gpu.h2d(dx, y)
        gpu.graph_launch(graph)
        got = gpu.download(dq, np.float32, (n, H, hd))
        calls()
        np.testing.assert_array_equal(gpu.download(dq, np.float32, (n, H, hd)), got)
        c.k[:], c.v[:], c.ks[:], c.vs[:] = c.pull()
        pos = np.arange(at, at + n)
        q = ref.rotate(y[:, :D].reshape(-1, H, hd), tab[pos], hd, 1)
        rows = [0, 1, 45, n - 1]
        K, V = c.values()
        close(got[rows], np.stack([ref.attend(q[i], K, V, 1, at + i + 1, 0.09) for i in rows]))
    gpu.graph_destroy(graph)
    for b in bufs:
        b.free()
    c.free()


def _dummy(gpu, c):
    return c.bufs[0], 128, c.bufs[1], 128


# ── together ──

def test_conversation(gpu):
    """Prompts of three sequences appended and attended, then tokens one by one, as a forward makes the calls; every
    output against float64 over the keys and values that the cache stands for, and the cache against the fp32 rows."""
    hd, kvh, H, max_seq = 128, 2, 14, 150
    D, KV = H * hd, kvh * hd
    rng = np.random.default_rng(20)
    scale, tab = 1 / math.sqrt(hd), ref.table(max_seq, hd)
    dt = gpu.upload(tab)
    rope = Rope(dt.ptr, max_seq, hd, 0)
    for kind in KINDS:
        c = ref.Cache(gpu, kind, 4, max_seq, kvh, hd, fill=0)
        lens, slot = [33, 1, 100], np.array([3, 0, 2], np.int32)
        n = sum(lens)
        tok_slot, tok_pos = np.repeat(slot, lens), np.concatenate([np.arange(m) for m in lens]).astype(np.int32)
        x = rng.standard_normal((n, D + 2 * KV)).astype(np.float32)
        bufs = [gpu.upload(x), i32(gpu, tok_slot), i32(gpu, tok_pos), gpu.alloc(4 * n * D), gpu.alloc(4 * n * D)]
        dx, ds, dp, dq, do = bufs

        def append(x, slot, pos):
            k = ref.rotate(x[:, D:D + KV].reshape(-1, kvh, hd), tab[pos], hd, 0)
            c.k[slot, :, pos], c.ks[slot, :, pos] = ref.rows(k, kind)
            c.v[slot, :, pos], c.vs[slot, :, pos] = ref.rows(x[:, D + KV:].reshape(-1, kvh, hd), kind)
            return ref.rotate(x[:, :D].reshape(-1, H, hd), tab[pos], hd, 0)

        ld = D + 2 * KV
        gpu.kv_append(c.kv, ds, dp, n, dx.offset(4 * D), dx.offset(4 * (D + KV)), ld, rope, dx, dq, H, ld, D)
        host = [np.array(a, np.int32) for a in (slot, [0, 0, 0], lens)]
        gpu.attn_prompt(do, D, dq, D, c.kv, *host, 3, H, scale)
        q = append(x, tok_slot, tok_pos)
        close(gpu.download(do, np.float32, (n, H, hd)), want_prompt(c, q, slot, [0, 0, 0], lens, scale))
        dl = i32(gpu, [0, 0, 0])
        for step in range(3):
            pos = np.array([m + step for m in lens], np.int32)
            y = rng.standard_normal((3, ld)).astype(np.float32)
            gpu.h2d(dx, y)
            gpu.h2d(ds, slot)
            gpu.h2d(dp, pos)
            gpu.h2d(dl, pos + 1)
            gpu.kv_append(c.kv, ds, dp, 3, dx.offset(4 * D), dx.offset(4 * (D + KV)), ld, rope, dx, dq, H, ld, D)
            gpu.attn_decode(do, D, dq, D, c.kv, ds, dl, 3, H, scale)
            q = append(y, slot, pos)
            close(gpu.download(do, np.float32, (3, H, hd)), want_decode(c, q, slot, pos + 1, scale))
        for b in bufs + [dl]:
            b.free()
        c.free()
    dt.free()


@pytest.mark.parametrize("kind", KINDS)
def test_captured(gpu, kind):
    """A step captured and replayed follows the device's slots, positions and lengths, with eager work in between."""
    hd, kvh, H, max_seq, n = 128, 2, 14, 700, 5
    D, KV = H * hd, kvh * hd
    ld = D + 2 * KV
    rng = np.random.default_rng(30)
    c = ref.Cache(gpu, kind, n + 1, max_seq, kvh, hd, rng)
    tab = ref.table(max_seq, hd)
    x = rng.standard_normal((n, ld)).astype(np.float32)
    bufs = [gpu.upload(x), i32(gpu, range(n)), i32(gpu, [0] * n), i32(gpu, [0] * n), gpu.alloc(4 * n * D),
            gpu.alloc(4 * n * D), gpu.upload(tab)]
    dx, ds, dp, dl, dq, do, dt = bufs
    rope = Rope(dt.ptr, max_seq, hd, 0)

    def step():
        gpu.kv_append(c.kv, ds, dp, n, dx.offset(4 * D), dx.offset(4 * (D + KV)), ld, rope, dx, dq, H, ld, D)
        gpu.attn_decode(do, D, dq, D, c.kv, ds, dl, n, H, 0.09, n, 64)

    step()   # the workspaces exist before the capture
    gpu.capture_begin()
    step()
    graph = gpu.capture_end()
    for r in range(4):
        pos = np.array([100 + r, 690 + r, 64, 300 - r, 65 + r], np.int32)
        slot = np.roll(np.arange(n, dtype=np.int32), r)
        y = rng.standard_normal((n, ld)).astype(np.float32)
        for b, a in ((dx, y), (ds, slot), (dp, pos), (dl, pos + 1)):
            gpu.h2d(b, a)
        gpu.graph_launch(graph)
        got = gpu.download(do, np.float32, (n, H, hd))
        step()
        np.testing.assert_array_equal(gpu.download(do, np.float32, (n, H, hd)), got)
        k = ref.rotate(y[:, D:D + KV].reshape(-1, kvh, hd), tab[pos], hd, 0)
        c.k[:], c.v[:], c.ks[:], c.vs[:] = c.pull()
        q = ref.rotate(y[:, :D].reshape(-1, H, hd), tab[pos], hd, 0)
        np.testing.assert_array_equal(c.k[slot, :, pos], ref.rows(k, kind)[0])
        close(got, want_decode(c, q, slot, pos + 1, 0.09, n, 64))
    gpu.graph_destroy(graph)
    for b in bufs:
        b.free()
    c.free()


def test_calls_repeat_themselves(gpu):
    """The same call, the same bits, whatever ran before it."""
    rng = np.random.default_rng(40)
    c = ref.Cache(gpu, KV_Q8, 9, 3000, 4, 128, rng)
    lens = [3000, 17, 2500, 64, 1, 2999, 1000, 1500]
    q = rng.standard_normal((8, 28, 128)).astype(np.float32)
    first = run_decode(gpu, c, q, None, lens, 0.09, 8, 900)
    qp = rng.standard_normal((300, 28, 128)).astype(np.float32)
    p1 = run_prompt(gpu, c, qp, None, [0, 2000], [100, 200], 0.09)
    np.testing.assert_array_equal(run_decode(gpu, c, q, None, lens, 0.09, 8, 900), first)
    np.testing.assert_array_equal(run_prompt(gpu, c, qp, None, [0, 2000], [100, 200], 0.09), p1)
    c.free()


def test_refused_calls_say_why(gpu):
    c = ref.Cache(gpu, KV_Q8, 2, 64, 1, 64, fill=0)
    with pytest.raises(HakoGpuError, match="query heads"):
        gpu.attn_decode(c.bufs[0], 1088, c.bufs[0], 1088, c.kv, None, c.bufs[2], 1, 17, 1.0)
    with pytest.raises(HakoGpuError, match="positions"):
        gpu.attn_prompt(c.bufs[0], 64, c.bufs[1], 64, c.kv, None, np.array([60], np.int32), np.array([5], np.int32), 1, 1, 1.0)
    c.free()


@pytest.mark.parametrize("kind", KINDS)
def test_two_graphs_and_a_growing_workspace(gpu, kind):
    """A captured call, a call that needs a larger workspace, a second captured one, and replays of both in turn, with eager
    calls and a read-back captured too: each answers as the eager call on the same inputs."""
    rng = np.random.default_rng(70)
    small = ref.Cache(gpu, kind, 3, 900, 2, 64, rng)
    large = ref.Cache(gpu, kind, 1, 131072 if kind == KV_Q8 else 140000, 4, 64, fill=0)
    n, H, m = 3, 8, 128
    lens = [900, 333, 1]
    dq, do, dl = gpu.alloc(4 * n * H * 64), gpu.alloc(4 * n * H * 64), i32(gpu, lens)
    ds, dp, dk = i32(gpu, [0, 1, 2]), i32(gpu, [5, 332, 0]), gpu.alloc(4 * n * 2 * 64)
    bq, bo, bl, bs = gpu.upload(rng.standard_normal((m, 64, 64)).astype(np.float32)), gpu.alloc(4 * m * 64 * 64), i32(gpu, [40] * m), i32(gpu, [0] * m)
    q = rng.standard_normal((n, H, 64)).astype(np.float32)

    def one():
        gpu.attn_decode(do, H * 64, dq, H * 64, small.kv, None, dl, n, H, 0.125)

    def two():
        gpu.attn_decode(do, H * 64, dq, H * 64, small.kv, None, dl, n, H, 0.125, 2, 100)
        gpu.kv_read(small.kv, ds, dp, n, dk, None, 2 * 64)

    def captured(call):
        call()
        gpu.capture_begin()
        call()
        return gpu.capture_end()

    def of(x):
        return gpu.download(x, np.float32, (n, H if x is do else 2, 64))

    gpu.h2d(dq, q)
    first = captured(one)
    gpu.attn_decode(bo, 64 * 64, bq, 64 * 64, large.kv, bs, bl, m, 64, 0.125)   # 64 records a head
    second = captured(two)
    for r in range(3):
        q = rng.standard_normal((n, H, 64)).astype(np.float32)
        gpu.h2d(dq, q)
        gpu.graph_launch(first)
        got = of(do)
        close(got, want_decode(small, q, None, lens, 0.125))
        gpu.graph_launch(second)
        got2, rows = of(do), of(dk)
        close(got2, want_decode(small, q, None, lens, 0.125, 2, 100))
        np.testing.assert_array_equal(rows, np.stack([small.k[s, :, p].astype(np.float32) * small.ks[s, :, p, None] for s, p in ((0, 5), (1, 332), (2, 0))]))
        one()
        np.testing.assert_array_equal(of(do), got)
        two()
        np.testing.assert_array_equal(of(do), got2)
    for g in (first, second):
        gpu.graph_destroy(g)
    for b in (dq, do, dl, ds, dp, dk, bq, bo, bl, bs):
        b.free()
    small.free()
    large.free()
