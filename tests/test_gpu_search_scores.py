"""Windows and drafted trees over keys and values of any size: the inputs, bound and derivation of
test_gpu_attn_scores.py's ties. One key beats all others by a wide margin at many positions, its scores round nowhere,
and a row's answer is the mean of the value rows at those of these positions that it sees."""
import numpy as np
import pytest

from hako_amd.gpu import KV_F16, KV_Q8
from test_gpu_attn_scores import TIES, dominated, rows_close, unit_scale
from test_gpu_tree import ancestors, masks, random_tree, run_tree
from test_gpu_window import run_decode, run_prompt

pytestmark = pytest.mark.gpu

TUNE_ATTN_PROMPT = 21
KINDS = [KV_Q8, KV_F16]
AT = [0, 5, 31, 32, 63, 64, 100, 127, 129, 200, 255, 256, 300, 511, 640, 900, 1023, 1024, 1100]


def mean_at(c, slot, positions, G):
    """positions: those that a row sees."""
    at = [p for p in AT if p in positions]
    return np.repeat(c.V[slot][:, at].mean(1), G, 0)


def in_sight(t, window, sinks):
    return {p for p in range(t + 1) if p > t - window or p < sinks}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", TIES, ids=str)
@pytest.mark.parametrize("flip", [False, True], ids=["large", "negative"])
def test_window_ties(gpu, kind, size, flip):
    scale = -unit_scale() if flip else unit_scale()
    c, q = dominated(gpu, kind, 5, 1200, 1, 64, size, AT, flip)
    lens = [1200, 1, 40, 700, 1101]
    for window, sinks in ((130, 3), (800, 70)):
        want = np.stack([mean_at(c, s, in_sight(m - 1, window, sinks), 4) for s, m in enumerate(lens)])
        rows_close(run_decode(gpu, c, q[:5], None, lens, scale, window, sinks), want)
    start, n = [0, 1000, 60], [100, 130, 70]
    for knob in (1, 2, 3):
        gpu.tune(TUNE_ATTN_PROMPT, knob)
        for window, sinks in ((90, 3), (500, 70)):
            want = [mean_at(c, s, in_sight(a + i, window, sinks), 4) for s, (a, m) in enumerate(zip(start, n)) for i in range(m)]
            rows_close(run_prompt(gpu, c, q, None, start, n, scale, window, sinks), np.stack(want))
    gpu.tune(TUNE_ATTN_PROMPT, 0)
    c.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", TIES, ids=str)
@pytest.mark.parametrize("flip", [False, True], ids=["large", "negative"])
def test_tree_ties(gpu, kind, size, flip):
    """Many parts and few (both joins), winners among the text's and the tree's rows."""
    scale = -unit_scale() if flip else unit_scale()
    c, q = dominated(gpu, kind, 5, 1200, 1, 128, size, AT, flip)
    rng = np.random.default_rng(6)
    for base, N in (([1018], 20), ([1018, 250, 1, 60, 1160], 30)):
        sets = [ancestors(random_tree(rng, N, N)) for _ in base]
        want = [mean_at(c, s, set(range(b)) | {b + i for i in sets[s][j]}, 4) for s, b in enumerate(base) for j in range(N)]
        for knob in (1, 2, 3):
            gpu.tune(TUNE_ATTN_PROMPT, knob)
            got = run_tree(gpu, c, q[:len(base) * N], None, base, np.stack([masks(s) for s in sets]), N, scale)
            rows_close(got.reshape(len(want), *q.shape[1:]), np.stack(want))
    gpu.tune(TUNE_ATTN_PROMPT, 0)
    c.free()
