"""Attention over keys and values of any size in 2^-80..2^80: scores of any size a float holds, value rows of any size.

Two kinds of inputs, every kernel (single tokens in one part and in several,
over a shared prefix, prompts by the direct and the tiled kernel):

* One key row that beats all others by a wide margin for every query, at many
  positions, so that the same score comes up in different steps, waves, parts
  and kernels. Queries of 1, 2 and 3, codes of one size and a scale that makes
  scale * log2(e) a power of two leave nothing to round in those scores, in any
  order of the sum, so the answer is the mean of the value rows at those
  positions the token sees, whatever the scores' size: 1e-5 of the row's largest
  output, as everywhere else.

* N(0, 1) queries and keys times a power of two. A score of head_dim products
  carries an error: 2^-22 of each product (the query's two halves), and 2^-24
  of the partial sums in 2 * head_dim / 16 steps of the matrix cores, so at
  most 2^-22 + 16 * 2^-24 of sum |q_d k_d|, with the two roundings of its
  factors below 2^-19 of it: d. Then a weight is off by a factor of at most
  exp(2 d) either way and not above 1, and an output by the sum over p of what
  that makes of |w_p|, times |v_p|; 1e-5 of the row's largest output on top.
  Where the two largest scores lie closer than d, that allows any mix of the
  two; where they do not, it asks for the right row.
"""
import numpy as np
import pytest

import attn_ref as ref
from hako_amd.gpu import KV_F16, KV_Q8
from test_gpu_attn import prompt_kernel, run_decode, run_prompt   # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

KINDS = [KV_Q8, KV_F16]
SIZES = [(0, 17), (10, 17), (16, 30), (17, 60), (19, -50), (22, 3), (24, 40), (26, 0), (30, 17), (40, 30), (60, 60),
         (60, -50), (72, 70), (-60, 60)]
TIES = [s for s in SIZES if s[0] >= 10]   # (there the others' weights are below e^-10000)


def unit_scale():
    """A float32 whose product with float32 log2(e) rounds to 1/8."""
    s = np.float32(0.125 / np.log2(np.e))
    for _ in range(4):
        s = np.nextafter(s, np.float32(0))
    while np.float32(s * np.float32(np.log2(np.e))) < np.float32(0.125):
        s = np.nextafter(s, np.float32(1))
    assert np.float32(s * np.float32(np.log2(np.e))) == np.float32(0.125)
    return float(s)


def rows_close(got, want, more=0.0):
    assert np.isfinite(got).all()
    off = np.abs(got - want) - 1e-5 * np.abs(want).max(-1, keepdims=True) - more
    assert (off <= 0).all(), f"{(off > 0).any(-1).sum()} rows, up to {(np.abs(got - want) / np.abs(want).max(-1, keepdims=True)).max():.3g}"


def dominated(gpu, kind, slots, max_seq, kvh, hd, size, at, flip):
    """A cache whose rows at positions `at` are the winning key; value rows of several sizes, the largest 2^size[1]."""
    rng = np.random.default_rng(100 * size[0] + size[1])
    c = ref.Cache(gpu, kind, slots, max_seq, kvh, hd, rng)
    # every query is positive: keys of all 1 against keys below 1/4, or, with a negative scale, keys of 1/16 against ones
    # of 1/4 to 1
    x = rng.uniform(0.25, 1, c.k.shape) if flip else rng.uniform(-0.25, 0.25, c.k.shape)
    x[:, :, at] = 1 / 16 if flip else 1
    c.k, c.ks = ref.rows(np.ldexp(x, size[0]), kind)
    v = np.ldexp(rng.standard_normal(c.v.shape), size[1])
    c.v, c.vs = ref.rows(v * 2.0 ** -(np.arange(max_seq) // 37 % 4 * 9)[None, None, :, None], kind)
    c.push()
    c.V = c.values()[1]
    q = rng.integers(1, 4, (300, 4 * kvh, hd)).astype(np.float32)
    return c, q


def mean_of_seen(c, slot, end, at, G, ps=0, pl=0):
    V = c.V
    at = np.asarray(at)
    at = at[at < end]
    rows = np.where((at < pl)[:, None, None], V[ps][:, at].transpose(1, 0, 2), V[slot][:, at].transpose(1, 0, 2))
    return np.repeat(rows.mean(0), G, 0)


AT = [0, 5, 31, 32, 63, 64, 100, 127, 129, 200, 255, 256, 300, 511, 640, 900, 1023, 1024, 1100]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", TIES, ids=str)
@pytest.mark.parametrize("flip", [False, True], ids=["large", "negative"])
def test_decode_ties(gpu, kind, size, flip):
    c, q = dominated(gpu, kind, 6, 1200, 2, 128, size, AT, flip)
    scale = -unit_scale() if flip else unit_scale()
    lens = [1200, 1, 40, 700, 1101]
    want = np.stack([mean_of_seen(c, s, m, AT, 4) for s, m in enumerate(lens)])
    rows_close(run_decode(gpu, c, q[:5], None, lens, scale), want)
    # over a prefix
    want = np.stack([mean_of_seen(c, s, m, AT, 4, 5, 650) for s, m in enumerate(lens)])
    rows_close(run_decode(gpu, c, q[:5], None, lens, scale, 5, 650), want)
    # in one part, many sequences
    slot, lens = [i % 6 for i in range(300)], [1 + (i * 41) % 1200 for i in range(300)]
    want = np.stack([mean_of_seen(c, s, m, AT, 4) for s, m in zip(slot, lens)])
    rows_close(run_decode(gpu, c, q, slot, lens, scale), want)
    c.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", TIES, ids=str)
@pytest.mark.parametrize("flip", [False, True], ids=["large", "negative"])
def test_prompt_ties(gpu, prompt_kernel, kind, size, flip):   # noqa: F811
    c, q = dominated(gpu, kind, 4, 1200, 1, 64, size, AT, flip)
    scale = -unit_scale() if flip else unit_scale()
    start, lens = [0, 1000, 60], [100, 130, 70]
    for ps, pl in ((0, 0), (3, 77)):
        want = [mean_of_seen(c, s, a + i + 1, AT, 4, ps, pl) for s, (a, m) in enumerate(zip(start, lens)) for i in range(m)]
        rows_close(run_prompt(gpu, c, q, None, start, lens, scale, ps, pl), np.stack(want))
    c.free()


def bounded(c, q, slot, end, scale):
    """One token's output in float64, and how far scores' errors may move it."""
    K, V = (x[slot, :, :end] for x in c.values())
    H, hd = q.shape
    G = H // K.shape[0]
    out, more = np.zeros((2, H, hd))
    for h in range(H):
        k, v, qd = K[h // G], V[h // G], q[h].astype(np.float64)
        s = k @ qd * scale
        d = 2.0 ** -19 * scale * (np.abs(k) @ np.abs(qd)).max()
        w = np.exp(s - s.max())
        w /= w.sum()
        grown = np.exp(np.minimum(0, s - s.max() - np.log(np.exp(s - s.max()).sum()) + 2 * d))
        lost = w * -np.expm1(-2 * d)
        out[h], more[h] = w @ v, np.maximum(grown - w, lost) @ np.abs(v)
    return out, more


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", SIZES + [(77, 77), (77, -77), (-77, 77), (-77, -77)], ids=str)   # (N(0, 1) to the ends of the range)
def test_random_keys(gpu, prompt_kernel, kind, size):   # noqa: F811
    rng = np.random.default_rng(size[0] + 77)
    c = ref.Cache(gpu, kind, 3, 700, 2, 128, rng)
    c.ks *= np.float32(2.0 ** size[0])
    c.vs *= np.float32(2.0 ** size[1])
    c.push()
    q = rng.standard_normal((90, 6, 128)).astype(np.float32)
    lens = [700, 333, 64]
    if prompt_kernel == 0:
        want, more = zip(*(bounded(c, q[s], s, m, 0.09) for s, m in enumerate(lens)))
        rows_close(run_decode(gpu, c, q[:3], None, lens, 0.09), np.stack(want), np.stack(more))
    start, lens = [0, 600], [40, 50]
    want, more = zip(*(bounded(c, q[i], int(i >= 40), i + 1 if i < 40 else 560 + i + 1, 0.09) for i in range(90)))
    rows_close(run_prompt(gpu, c, q, None, start, lens, 0.09), np.stack(want), np.stack(more))
    c.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [30, 60])
def test_later_rows_do_not_count(gpu, prompt_kernel, kind, size):   # noqa: F811
    """Scores of a size that the other rows of a wave do not have: those rows' outputs do not move by a bit."""
    rng = np.random.default_rng(6)
    c = ref.Cache(gpu, kind, 2, 200, 1, 128, rng)
    start, lens, at = [0, 30], [100, 71], 60
    q = rng.standard_normal((171, 4, 128)).astype(np.float32)
    before = [i for i in range(171) if (i if i < 100 else i - 70) < at]
    first = run_prompt(gpu, c, q, None, start, lens, 0.09)
    c.ks[:, :, at:] *= np.float32(2.0 ** size)
    c.vs[:, :, at:] *= np.float32(2.0 ** size)
    c.push()
    got = run_prompt(gpu, c, q, None, start, lens, 0.09)
    np.testing.assert_array_equal(got[before], first[before])
    want, more = zip(*(bounded(c, q[i], int(i >= 100), i + 1 if i < 100 else i - 69, 0.09) for i in range(171)))
    rows_close(got, np.stack(want), np.stack(more))
    c.free()
