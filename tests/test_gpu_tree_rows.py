"""Rows of the cache that no node of a drafted tree sees: a padded tree's, which nobody wrote. Whatever they hold, outputs
are those of the rows that are seen (float64, bound and derivation of test_gpu_attn.py)."""
import math

import numpy as np
import pytest

import attn_ref as ref
from hako_amd.gpu import KV_F16, KV_Q8
from test_gpu_tree import ancestors, attend, close, kernel, masks, random_tree, run_tree   # noqa: F401

pytestmark = pytest.mark.gpu


def spoil(c, slot, row):
    """What memory may hold before its first use: any bits."""
    code = (127, -127) if c.kind == KV_Q8 else (np.nan, np.inf)
    c.k[slot, :, row], c.v[slot, :, row] = code if row % 2 else code[::-1]
    c.ks[slot, :, row], c.vs[slot, :, row] = ((np.nan, 1.0), (1.0, 1.0), (np.inf, np.nan), (3e38, 3e38))[row % 4]


@pytest.mark.parametrize("kind", [KV_F16, KV_Q8])
@pytest.mark.parametrize("H,KVH,hd", [(28, 4, 128), (4, 2, 64), (16, 1, 64)])
@pytest.mark.parametrize("N", [2, 20, 64])
def test_padded_trees_over_unwritten_rows(gpu, kernel, kind, H, KVH, hd, N):   # noqa: F811
    rng = np.random.default_rng(N + H)
    base, max_seq = [0, 1, 30, 33, 63, 64, 100, 700], 800
    n = len(base)
    c = ref.Cache(gpu, kind, n, max_seq, KVH, hd, rng)
    K, V = c.values()
    sets = [ancestors(random_tree(rng, int(rng.integers(1, N)), N)) for _ in base]
    for i, b in enumerate(base):
        used = set().union(*sets[i])
        for row in range(b, max_seq):
            if row - b not in used:
                spoil(c, i, row)
    c.push()
    q = rng.standard_normal((n * N, H, hd)).astype(np.float32)
    got = run_tree(gpu, c, q, None, base, np.stack([masks(s) for s in sets]), N, 1 / math.sqrt(hd))
    for i in range(n):
        close(got[i], np.array([attend(q[i * N + j], K, V, i, base[i], sets[i][j], max_seq, 1 / math.sqrt(hd)) for j in range(N)]))
    c.free()


@pytest.mark.parametrize("prefix", [0, 500])
def test_nodes_missing_among_others(gpu, kernel, prefix):   # noqa: F811
    """Masks with holes, in parts and over a prefix: rows past the last node's, first ones and ones between them."""
    H, KVH, hd, N, max_seq = 16, 2, 128, 64, 2200
    rng = np.random.default_rng(prefix)
    base = [2000, 1990, 2100]
    n = len(base)
    c = ref.Cache(gpu, KV_F16, n + 1, max_seq, KVH, hd, rng)
    K, V = c.values()
    there = [{0, 3, 4, 31, 32, 40}, {1, 2, 62, 63}, {5}]
    seen = [[{i for i in t if i <= j} if j in t else set() for j in range(N)] for t in there]
    for i, b in enumerate(base):
        for row in range(b, max_seq):
            if row - b not in there[i]:
                spoil(c, i, row)
    c.push()
    q = rng.standard_normal((n * N, H, hd)).astype(np.float32)
    got = run_tree(gpu, c, q, None, base, np.stack([masks(s) for s in seen]), N, 0.09, (n, prefix))
    for i in range(n):
        close(got[i], np.array([attend(q[i * N + j], K, V, i, base[i], seen[i][j], max_seq, 0.09, n, prefix) for j in range(N)]))
    c.free()
