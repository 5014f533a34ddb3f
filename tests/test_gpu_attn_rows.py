"""Attention row by row: each token's query head against its own largest output in float64.

In a long causal prompt the first tokens' outputs are a hundred times the last
ones', so a bound by the largest output of the call says little of the long
rows. Here a row (token, query head) of up to 10^4 positions may be 1e-5 of its
own largest output off, and one that sees nothing is zeros. What goes into that
bound, for N(0, 1) queries, keys and values and scores of up to about 4:

* a weight's own error, from its score: the query's 22 bits over head_dim
  products 7e-8, the 2 head_dim / 16 partial sums' roundings 3e-7, the fused
  multiply-add and the exponential 3e-7; together 5e-7, independent from key to
  key, so it moves an output by that part of sqrt(sum w^2 v^2), which is the
  output's own size;
* the sums over n positions: 2 n / 16 roundings of partial sums that grow to the
  output like a random walk, 2^-25 sqrt(n / 16) of it, 7e-7 at 10^4; the sum of
  the weights, n / 2 additions in a lane, 2^-25 sqrt(n / 6), 1.2e-6.

That is 2.5e-6 in the root mean square at 10^4 positions, 1.5e-6 below 10^3;
the largest of a row's 128 outputs errs 2.6 of them and is itself 2.6 of its
row's. 1e-5 is four times that. Weights or queries without their low halves err
by 2^-12 and more (test_the_bound_sees_a_missing_half).
"""
import math

import numpy as np
import pytest

import attn_ref as ref
from hako_amd.gpu import KV_F16, KV_Q8
from test_gpu_attn import prompt_kernel, run_decode, run_prompt, want_decode, want_prompt   # noqa: F401 (a fixture)

KINDS = [KV_Q8, KV_F16]
TOL = 1e-5


def off(got, want):
    """The largest error of the rows of want, as a part of the row's largest output; rows of zeros have none."""
    top = np.abs(want).max(-1)
    assert np.isfinite(got).all() and (got[top == 0] == 0).all()
    return (np.abs(got - want).max(-1)[top > 0] / top[top > 0]).max()


@pytest.mark.parametrize("n", [64, 1000, 8000])
@pytest.mark.parametrize("half", ["weights", "queries"])
def test_the_bound_sees_a_missing_half(n, half):
    rng = np.random.default_rng(n)
    q, k, v = rng.standard_normal((16, 128)), rng.standard_normal((n, 128)), rng.standard_normal((n, 128))
    s = q @ k.T / math.sqrt(128)
    w = np.exp(s - s.max(1, keepdims=True))
    l = w.sum(1, keepdims=True)
    want = w @ v / l
    if half == "weights":
        got = w.astype(np.float16).astype(np.float64) @ v / l
    else:
        s = q.astype(np.float16).astype(np.float64) @ k.T / math.sqrt(128)
        w = np.exp(s - s.max(1, keepdims=True))
        got = w @ v / w.sum(1, keepdims=True)
    assert (np.abs(got - want).max(1) / np.abs(want).max(1)).min() > 3 * TOL


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,kvh,G,max_seq,lens,ps,pl", [
    (128, 2, 8, 9000, [9000, 1, 0, 33, 5000, 700], 0, 0), (128, 4, 7, 5000, [5000, 4097, 64, 1], 3, 3000),
    (64, 1, 16, 9999, [9999, 100], 1, 90), (128, 1, 1, 257, [257, 256, 0, 1], 0, 0)])
def test_decode(gpu, kind, hd, kvh, G, max_seq, lens, ps, pl):
    rng = np.random.default_rng(max_seq + hd)
    c = ref.Cache(gpu, kind, len(lens), max_seq, kvh, hd, rng)
    q = rng.standard_normal((len(lens), kvh * G, hd)).astype(np.float32)
    scale = 1 / math.sqrt(hd)
    assert off(run_decode(gpu, c, q, None, lens, scale, ps, pl), want_decode(c, q, None, lens, scale, ps, pl)) < TOL
    c.free()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,kvh,G,start,lens,prefix", [
    (128, 4, 7, [0, 500], [4500, 700], 0), (64, 1, 16, [0], [8100], 0), (128, 8, 4, [1000, 1000, 1000], [1500, 40, 900], 1000),
    (128, 2, 3, [0, 3000], [77, 200], 0), (64, 2, 5, [1, 8000], [130, 64], 40)])
def test_prompt(gpu, prompt_kernel, kind, hd, kvh, G, start, lens, prefix):   # noqa: F811
    if prompt_kernel == 1 and sum(lens) > 5000:
        pytest.skip("the tiled kernel's range")
    rng = np.random.default_rng(hd * G)
    n_seq, scale = len(lens), 1 / math.sqrt(hd)
    c = ref.Cache(gpu, kind, n_seq + 1, max(a + m for a, m in zip(start, lens)), kvh, hd, rng)
    q = rng.standard_normal((sum(lens), kvh * G, hd)).astype(np.float32)
    got = run_prompt(gpu, c, q, None, start, lens, scale, n_seq, prefix)
    K, V = c.values()
    row, at, want = 0, [], []
    for s, (a, m) in enumerate(zip(start, lens)):
        for i in {*range(0, m, max(1, m // 40)), min(1, m - 1), m - 1}:
            at.append(row + i)
            want.append(ref.attend(q[row + i], K, V, s, a + i + 1, scale, n_seq, prefix))
        row += m
    assert off(got[at], np.stack(want)) < TOL
    c.free()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [70, 20, -20, -70])
@pytest.mark.parametrize("first", [-9, -40, 9])
def test_values_of_two_sizes(gpu, prompt_kernel, kind, size, first):   # noqa: F811
    """Value rows before position 70 are 2^first of those after it: a row that sees the former alone is as exact as one
    that sees both."""
    rng = np.random.default_rng(size + 100)
    c = ref.Cache(gpu, kind, 1, 300, 2, 64, rng)
    c.vs *= np.float32(2.0 ** size)
    c.vs[:, :, :70] *= np.float32(2.0 ** (first if size > -70 else abs(first)))
    c.push()
    q = rng.standard_normal((90, 6, 64)).astype(np.float32)
    for start in (0, 45, 210):
        assert off(run_prompt(gpu, c, q, None, [start], [90], 0.125), want_prompt(c, q, None, [start], [90], 0.125)) < TOL
    for n in (40, 71, 300):
        assert off(run_decode(gpu, c, q[:1], None, [n], 0.125), want_decode(c, q[:1], None, [n], 0.125)) < TOL
    c.free()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_rows_that_see_nothing(gpu, kind):
    """Exact zeros in every path: one part, several, over a prefix, in place."""
    rng = np.random.default_rng(4)
    c = ref.Cache(gpu, kind, 6, 3000, 2, 128, rng)
    slot, lens = [0, 1, 2, 9, 4, -1], [3000, 0, -7, 100, 1, 5]
    q = rng.standard_normal((6, 14, 128)).astype(np.float32)
    for ps, pl, in_place in ((0, 0, False), (5, 500, False), (5, 500, True), (5, 3000, False)):
        want = want_decode(c, q, slot, lens, 0.09, ps, pl)
        assert (want[[1, 2, 3, 5]] == 0).all() and (want[[0, 4]] != 0).any((1, 2)).all()
        assert off(run_decode(gpu, c, q, slot, lens, 0.09, ps, pl, pad=4, in_place=in_place), want) < TOL
    c.free()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_queries_that_are_not_finite(gpu, prompt_kernel, kind):   # noqa: F811
    """A query head with a NaN or an infinity answers NaN; the other heads and tokens do not move by a bit."""
    rng = np.random.default_rng(8)
    c = ref.Cache(gpu, kind, 3, 900, 2, 128, rng)
    q = rng.standard_normal((150, 8, 128)).astype(np.float32)
    bad = [(0, 0, np.nan), (1, 3, np.inf), (2, 7, -np.inf), (100, 5, np.nan), (149, 0, np.inf)]
    hurt = q.copy()
    for t, h, x in bad:
        hurt[t, h, (t + h) % 128] = x
    where = np.zeros(q.shape[:2], bool)
    for t, h, _ in bad:
        where[t, h] = True

    def check(first, got):
        assert np.isnan(got[where[:len(got)]]).all()
        np.testing.assert_array_equal(got[~where[:len(got)]], first[~where[:len(got)]])
        assert np.isfinite(first).all()

    for ps, pl in ((0, 0), (2, 300)):
        check(*(run_prompt(gpu, c, x, None, [0, 700], [70, 80], 0.09, ps, pl) for x in (q, hurt)))
        check(*(run_decode(gpu, c, x[:3], None, [900, 400, 30], 0.09, ps, pl) for x in (q, hurt)))
    c.free()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale", [-0.09, 0.0])
def test_scales(gpu, prompt_kernel, kind, scale):   # noqa: F811
    """A negative scale, and 0: the mean of the values seen."""
    rng = np.random.default_rng(9)
    c = ref.Cache(gpu, kind, 2, 500, 2, 64, rng)
    q = rng.standard_normal((130, 6, 64)).astype(np.float32)
    assert off(run_prompt(gpu, c, q, None, [0, 440], [70, 60], scale), want_prompt(c, q, None, [0, 440], [70, 60], scale)) < TOL
    assert off(run_decode(gpu, c, q[:2], None, [500, 3], scale), want_decode(c, q[:2], None, [500, 3], scale)) < TOL
    c.free()


@pytest.mark.gpu
def test_many_prompts_in_place(gpu, prompt_kernel):   # noqa: F811
    """More sequences than a launch takes, in place, over a prefix: a launch does not touch the rows of the others."""
    rng = np.random.default_rng(10)
    n = 130
    c = ref.Cache(gpu, KV_F16, 11, 400, 1, 64, rng)
    lens, start = [1 + (i * 7) % 23 for i in range(n)], [(i * 31) % 370 for i in range(n)]
    slot = [i % 10 for i in range(n)]
    q = rng.standard_normal((sum(lens), 4, 64)).astype(np.float32)
    want = want_prompt(c, q, slot, start, lens, 0.125, 10, 150)
    assert off(run_prompt(gpu, c, q, slot, start, lens, 0.125, 10, 150, pad=4, in_place=True), want) < TOL
    c.free()
